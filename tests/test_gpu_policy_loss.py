"""The clipped policy loss and its gradient against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
import vocabulary_reference as V
from minml_amd import core as ml
from test_gpu_gated import check_guards, guarded

pytestmark = pytest.mark.gpu
CLIP, KL_WEIGHT, CLASSES = (0.2, 0.28), float(np.float32(0.04)), 1000


def inputs(rng, sequences, length, per_token=False):
    old = rng.exponential(1.0, (sequences, length)).astype(np.float32)
    nll = np.maximum(old + rng.normal(0, 0.3, old.shape), 0).astype(np.float32)
    reference = np.maximum(old + rng.normal(0, 0.6, old.shape), 0).astype(np.float32)
    advantages = rng.standard_normal((sequences, length) if per_token else sequences).astype(np.float32)
    targets = rng.integers(0, CLASSES, old.shape)
    places = np.arange(length)[None]
    begin = (rng.random((sequences, 1)) * 0.3 * length).astype(int)
    targets[(places < begin) | (places >= begin + (rng.random((sequences, 1)) * 1.2 * (length + 1)).astype(int))] = -1
    other = rng.random(old.shape) < 0.02
    targets[other] = rng.choice([-100, CLASSES, 2 ** 31 - 1, -2 ** 31], int(other.sum()))
    return nll, old, reference, advantages, targets.astype(np.int32)


class Loss:
    """The two calls with everything around them."""

    def __init__(self, ctx, nll, old, reference, advantages, targets, clip=CLIP, kl_weight=KL_WEIGHT, average="tokens"):
        self.ctx, self.clip, self.kl_weight = ctx, clip, kl_weight
        self.inputs = [None if a is None else guarded(ctx, a, "float32", np.nan) for a in (nll, old, reference, advantages)] + [ml.toDevice(ctx, targets)]
        sequences = nll.shape[0] if nll.ndim == 2 else 1
        self.loss, self.weights = (guarded(ctx, np.full(n, np.nan, np.float32), "float32", 9.0) for n in (4, sequences))
        space = V.workspace(ctx, ml.policyLossGetWorkspaceSize(ctx, self.inputs[0]))
        ml.policyLossForward(ctx, *self.inputs, CLASSES, clip, kl_weight, average, self.loss, self.weights, space)
        V.check_workspace(ctx, space)

    def gradient(self, dloss=None, beta=0.0, before=None):
        shape = self.inputs[0].shape
        dnll = guarded(self.ctx, np.full(shape, np.nan, np.float32) if before is None else before, "float32", 9.0)
        ml.policyLossBackward(self.ctx, *self.inputs, CLASSES, self.clip, self.kl_weight, self.weights, None if dloss is None else ml.toDevice(self.ctx, np.array([dloss], np.float32)), beta, dnll)
        check_guards(self.ctx, dnll, 9.0)
        return dnll.copyToHost(self.ctx)


def exact(nll, old, reference, advantages, targets, average, clip=CLIP, kl_weight=KL_WEIGHT):
    wide = lambda a: None if a is None else a.astype(np.float64)
    return V.policy(wide(nll), wide(old), wide(reference), wide(advantages), targets, CLASSES, clip, kl_weight, average)


# every way through: sequences by 8 threads, a wavefront, a workgroup, in chunks; tokens one by one and in fours; several sequences to a workgroup, more than the groups
SIZES = [(1, 1), (3, 2), (1, 3), (2, 4), (40, 5), (9000, 3), (5000, 7), (33, 64), (7, 65), (300, 113), (4, 1024), (3000, 40), (5, 1025), (600, 1030), (2, 8191), (1, 8192), (3, 20001), (1, 300001)]


@pytest.mark.parametrize("average", ["tokens", "sequences"])
@pytest.mark.parametrize("sequences,length", SIZES)
def test_loss_and_gradient(ctx, sequences, length, average):
    rng = np.random.default_rng(sequences * 10007 + length)
    for per_token, with_reference in ((False, True), (True, True), (True, False)):
        data = list(inputs(rng, sequences, length, per_token))
        if not with_reference:
            data[2] = None
        step = Loss(ctx, *data, average=average)
        (loss, weights, gradient), (loss_off, weights_off, gradient_off) = exact(*data, average)
        assert R.worst(step.loss.copyToHost(ctx), loss, loss_off) <= 1
        assert R.worst(step.weights.copyToHost(ctx), weights, weights_off + 1e-300) <= 1
        check_guards(ctx, step.loss, 9.0)
        check_guards(ctx, step.weights, 9.0)
        assert R.worst(step.gradient(), gradient, gradient_off) <= 1
        before = rng.standard_normal(gradient.shape).astype(np.float32)
        assert R.worst(step.gradient(512.0, -0.5, before), 512 * gradient - 0.5 * before, 512 * gradient_off + 2 * R.rounded(before, "float32")) <= 1


def test_one_sequence_without_leading_dimension(ctx):
    rng = np.random.default_rng(1)
    data = inputs(rng, 1, 70)
    both = [Loss(ctx, *data), Loss(ctx, *(a.reshape(-1) for a in data))]
    assert np.array_equal(both[0].loss.copyToHost(ctx), both[1].loss.copyToHost(ctx))
    assert np.array_equal(both[0].gradient()[0], both[1].gradient())


@pytest.mark.parametrize("average", ["tokens", "sequences"])
def test_what_masked_tokens_hold_reaches_nothing(ctx, average):
    rng = np.random.default_rng(2)
    for sequences, length in ((5, 3), (40, 90), (3, 9000)):
        for per_token in (False, True):
            data = list(inputs(rng, sequences, length, per_token))
            data[4][1] = -1  # a sequence without any token
            masked = (data[4] < 0) | (data[4] >= CLASSES)
            clean = Loss(ctx, *data, average=average)
            for i in (0, 1, 2) + ((3,) if per_token else ()):
                data[i] = np.where(masked, rng.choice([np.nan, np.inf, -np.inf, 1e38], data[i].shape), data[i]).astype(np.float32)
            if not per_token:
                data[3][1] = np.nan
            dirty = Loss(ctx, *data, average=average)
            assert np.array_equal(clean.loss.copyToHost(ctx), dirty.loss.copyToHost(ctx)) and np.array_equal(clean.weights.copyToHost(ctx), dirty.weights.copyToHost(ctx))
            assert np.isfinite(clean.loss.copyToHost(ctx)).all() and clean.weights.copyToHost(ctx)[1] == 0
            gradient = dirty.gradient()
            assert np.array_equal(gradient, clean.gradient()) and (gradient[masked] == 0).all()


@pytest.mark.parametrize("average", ["tokens", "sequences"])
def test_no_tokens_at_all(ctx, average):
    for shape in ((3, 50), (2, 2), (4, 0), (0, 7), (1, 10000)):
        data = [np.ones(shape, np.float32)] * 3 + [np.ones(shape[0], np.float32), np.full(shape, -1, np.int32)]
        step = Loss(ctx, *data, average=average)
        assert (step.loss.copyToHost(ctx) == 0).all() and (step.weights.copyToHost(ctx) == 0).all() and (step.gradient() == 0).all()


def test_tokens_at_the_border_of_the_clip(ctx):
    """Neighbouring numbers on both sides of the border, for either sign of the advantage; an advantage of 0; a clip of 0 at equal likelihoods; a lower border that nothing reaches; no upper border."""
    for clip in ((0.2, 0.28), (0.0, 0.0), (1.0, np.inf), (1.5, 0.1)):
        old = np.float32(4.0) + np.zeros((6, 64), np.float32)
        with np.errstate(divide="ignore"):
            at = [np.log1p(clip[1]), np.log1p(-clip[0]) if clip[0] < 1 else -30.0]
        nll = old.copy()
        for row, border in ((0, at[0]), (1, at[0]), (2, at[1]), (3, at[1])):
            if np.isfinite(border):
                middle = np.float32(4.0 - border)
                nll[row] = middle + np.arange(-32, 32) * np.spacing(middle)
        advantages = np.array([1, -1, 1, -1, 0, 1], np.float32)
        targets = np.zeros(old.shape, np.int32)
        step = Loss(ctx, nll, old, None, advantages, targets, clip=clip)
        (loss, _, gradient), (loss_off, _, gradient_off) = exact(nll, old, None, advantages, targets, "tokens", clip=clip)
        got = step.gradient()
        assert np.array_equal(got == 0, gradient == 0)
        assert R.worst(got, gradient, gradient_off) <= 1 and R.worst(step.loss.copyToHost(ctx), loss, loss_off) <= 1


def test_gradient_against_differences(ctx):
    """The gradient of the definition itself, away from the borders, by central differences in 64 bits."""
    rng = np.random.default_rng(3)
    data = [a.astype(np.float64) if a.dtype == np.float32 else a for a in inputs(rng, 2, 9, True)]
    gradient = exact(*data, "sequences")[0][2]
    for s in range(2):
        for t in range(9):
            d = data[1][s, t] - data[0][s, t]
            if min(abs(d - np.log1p(CLIP[1])), abs(d - np.log1p(-CLIP[0]))) < 1e-4:
                continue
            values = []
            for step in (1e-5, -1e-5):
                nll = data[0].copy()
                nll[s, t] += step
                values.append(exact(nll, *data[1:], "sequences")[0][0][0])
            assert abs((values[0] - values[1]) / 2e-5 - gradient[s, t]) < 1e-8


def test_tensors_that_begin_at_any_element(ctx):
    rng = np.random.default_rng(4)
    for sequences, length in ((3, 61), (300, 77), (2, 9001)):
        data = inputs(rng, sequences, length, True)
        plain = Loss(ctx, *data)
        shifted = [ml.toDevice(ctx, np.concatenate([a.reshape(-1)[:1], a.reshape(-1)])).view(a.shape, 1) for a in data]
        loss, weights, dnll = ml.Tensor((5,), "float32").view((4,), 1), ml.Tensor((sequences + 1,), "float32").view((sequences,), 1), ml.Tensor((sequences * length + 1,), "float32").view((sequences, length), 1)
        space = ml.Tensor((max(1, ml.policyLossGetWorkspaceSize(ctx, shifted[0])),), "uint8")
        ml.policyLossForward(ctx, *shifted, CLASSES, CLIP, KL_WEIGHT, "tokens", loss, weights, space)
        ml.policyLossBackward(ctx, *shifted, CLASSES, CLIP, KL_WEIGHT, weights, None, 0.0, dnll)
        assert np.array_equal(loss.copyToHost(ctx), plain.loss.copyToHost(ctx)) and np.array_equal(weights.copyToHost(ctx), plain.weights.copyToHost(ctx))
        assert np.array_equal(dnll.copyToHost(ctx), plain.gradient())


def test_ratios_beyond_fp32(ctx):
    """exp(100) is no number of fp32: an advantage of 0 makes nothing of it, a positive one is held by the clip, a negative one counts with what the product is, if that is a number again; whole sequences, one after the other,
    by 8 threads, by a wavefront and by a workgroup."""
    advantages = np.array([0, 1, -2.0 ** -70, 0, 2, -2.0 ** -100], np.float32)
    for length in (3, 50, 500, 2000):
        for per_token in (False, True):
            old, nll = np.repeat(np.array([[101, 101, 101, 1, 1, 131], [1, 1, 1, 121, 121, 1]], np.float32)[:, :, None], length, 2)
            given = np.repeat(advantages[:, None], length, 1) if per_token else advantages
            targets = np.zeros(old.shape, np.int32)
            for average in ("tokens", "sequences"):
                step = Loss(ctx, nll, old, None, given, targets, average=average)
                loss, _, gradient = exact(nll, old, None, given, targets, average)[0]
                assert np.isfinite(gradient).all() and (gradient[[0, 1, 3]] == 0).all() and abs(gradient[2]).min() > 0
                # an exponent of up to 130, rounded, an exponential, a product and the means, all of one sign beside the few clipped ones; nothing where it is 0
                assert R.worst(step.loss.copyToHost(ctx), loss, 146 * R.FP32 * abs(loss) + 1e-300) <= 1 and R.worst(step.gradient(), gradient, 146 * R.FP32 * abs(gradient) + 2.0 ** -140) <= 1


def test_infinite_ratios_without_advantage(ctx):
    """A token that was impossible when it was sampled (old_nll inf) or is now (nll inf): nothing without an advantage, but a likelihood that is no number is none."""
    old, nll = np.array([[np.inf, 1, 1, 1]], np.float32), np.array([[1, np.inf, 1, 2]], np.float32)
    advantages, targets = np.zeros((1, 4), np.float32), np.zeros((1, 4), np.int32)
    step = Loss(ctx, nll, old, None, advantages, targets)
    assert (step.loss.copyToHost(ctx) == 0).all() and (step.gradient() == 0).all()
    nll[0, 2] = np.nan
    step = Loss(ctx, nll, old, None, advantages, targets)
    assert np.isnan(step.loss.copyToHost(ctx)[0]) and np.array_equal(np.isnan(step.gradient()), [[False, False, True, False]])


def test_divergences_beyond_fp32(ctx):
    """exp(q) - q - 1 of q = 100 is no number of fp32, but a small weight makes one of it; of an impossible token it is infinite, not undefined."""
    rng = np.random.default_rng(5)
    for length in (3, 50, 2000):
        nll = rng.uniform(0.5, 2, (4, length)).astype(np.float32)
        nll[1] += 100
        old, reference, advantages, targets = nll.copy(), np.ones(nll.shape, np.float32), np.ones(4, np.float32), np.zeros(nll.shape, np.int32)
        weight = float(np.float32(1e-20))
        step = Loss(ctx, nll, old, reference, advantages, targets, kl_weight=weight)
        (loss, _, gradient), (loss_off, _, gradient_off) = exact(nll, old, reference, advantages, targets, "tokens", kl_weight=weight)
        assert loss[0] > 1e20 and R.worst(step.gradient(), gradient, gradient_off) <= 1
        got = step.loss.copyToHost(ctx)
        assert got[2] == np.inf and R.worst(got[[0, 1, 3]], loss[[0, 1, 3]], loss_off[[0, 1, 3]]) <= 1
        nll[1, 0] = np.inf
        step = Loss(ctx, nll, old, reference, advantages, targets)
        assert np.array_equal(step.loss.copyToHost(ctx)[[0, 2]], [np.inf, np.inf])


@pytest.mark.parametrize("average", ["tokens", "sequences"])
def test_divergences_without_weight(ctx, average):
    """With a weight of 0 the reference has no part in the loss and its gradient, however far away it is: the bits are those of a call without one, and the mean divergence is given all the same."""
    rng = np.random.default_rng(6)
    for sequences, length in ((3, 3), (5, 60), (40, 700), (2, 9000)):
        data = list(inputs(rng, sequences, length))
        data[4][0, 0] = 1
        nothing = Loss(ctx, data[0], data[1], None, *data[3:], kl_weight=0.0, average=average)
        for far, mean in ((data[0] - 100, np.inf), (data[0] - 1000, np.inf), (np.full_like(data[0], -np.inf), np.inf), (np.full_like(data[0], np.nan), np.nan), (data[0] - 1, np.e - 2)):
            data[2] = far.astype(np.float32)
            step = Loss(ctx, *data, kl_weight=0.0, average=average)
            loss, want = step.loss.copyToHost(ctx), nothing.loss.copyToHost(ctx)
            assert np.array_equal(loss[[0, 1, 3]], want[[0, 1, 3]]) and np.isfinite(loss[0]) and np.array_equal(step.gradient(), nothing.gradient())
            # nll - 1 is rounded to fp32, by 2^-24 of numbers up to 8 beside a slope of e - 1
            assert (np.array_equal(loss[2], mean, equal_nan=True) if not np.isfinite(mean) else abs(loss[2] - mean) < 32 * R.FP32)
