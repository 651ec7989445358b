"""The operators as a training step uses them, one after the other: a block of a language or policy model of normalisation, gated dense layer, down projection and residual, then normalisation and the
cross entropy over many classes; and its gradients all the way back to the input."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml

pytestmark = pytest.mark.gpu
EPSILON = 1e-5


def parameters(rng, features, hidden, classes):
    return dict(w1=1 + 0.1 * rng.standard_normal(features), b1=0.1 * rng.standard_normal(features), wg=rng.standard_normal((2, hidden, features)) / np.sqrt(features),
                bg=0.1 * rng.standard_normal((2, hidden)), wd=rng.standard_normal((features, hidden)) / np.sqrt(hidden), w2=1 + 0.1 * rng.standard_normal(features),
                b2=0.1 * rng.standard_normal(features), wc=2 * rng.standard_normal((classes, features)) / np.sqrt(features), bc=0.1 * rng.standard_normal(classes))


class Step:
    """Everything a program keeps: tensors, workspaces, gradients. forward() and backward() are the calls it makes."""

    def __init__(self, ctx, x, targets, dloss, p, dtype):
        self.ctx = ctx
        rows, features = x.shape
        hidden, classes = p["wg"].shape[1], p["wc"].shape[0]
        dev = lambda a: ml.toDevice(ctx, R.bits(a, dtype))
        self.x, self.targets, self.dloss = dev(x), ml.toDevice(ctx, targets), ml.toDevice(ctx, dloss)
        self.p = {k: dev(v) for k, v in p.items()}
        new = lambda *s, d=dtype: ml.Tensor(s, d)
        self.n1, self.h, self.kept, self.res, self.n2 = new(rows, features), new(rows, hidden), new(rows, 2, hidden), new(rows, features), new(rows, features)
        self.loss, self.lse = new(rows, d="float32"), new(rows, d="float32")
        self.g = {k: new(*v.shape) for k, v in p.items()}
        self.dn2, self.dres, self.dh, self.dn1, self.dx = new(rows, features), new(rows, features), new(rows, hidden), new(rows, features), new(rows, features)
        size = max(ml.layerNormGetWorkspaceSize(ctx, self.x), ml.gatedDenseGetWorkspaceSize(ctx, self.n1, self.p["wg"], True), ml.gatedDenseGetWorkspaceSize(ctx, self.n1, self.p["wg"], False),
                   ml.linearCrossEntropyGetWorkspaceSize(ctx, self.n2, self.p["wc"], True))
        self.space = new(size, d="uint8")  # one workspace for all of them: the calls of a stream follow one another

    def forward(self):
        c, p = self.ctx, self.p
        ml.layerNormForward(c, self.x, p["w1"], p["b1"], self.n1, EPSILON)
        ml.gatedDenseForward(c, self.n1, p["wg"], p["bg"], self.h, self.kept, "silu", self.space)
        ml.gemm_ex(c, self.res, 1.0, "n", self.h, "t", p["wd"], 1.0, self.x, None, "linear")
        ml.layerNormForward(c, self.res, p["w2"], p["b2"], self.n2, EPSILON)
        ml.linearCrossEntropyForward(c, self.n2, p["wc"], p["bc"], self.targets, self.loss, self.lse, self.space)

    def backward(self):
        c, p, g = self.ctx, self.p, self.g
        ml.linearCrossEntropyBackward(c, self.n2, p["wc"], p["bc"], self.targets, self.lse, self.dloss, 0.0, self.dn2, 0.0, g["wc"], g["bc"], self.space)
        ml.layerNormBackward(c, self.res, p["w2"], self.dn2, 0.0, self.dres, 0.0, g["w2"], g["b2"], self.space, EPSILON)
        ml.gemm(c, "n", "n", self.dh, self.dres, p["wd"])
        ml.gemm(c, "t", "n", g["wd"], self.dres, self.h)
        ml.gatedDenseBackward(c, self.n1, p["wg"], self.kept, self.dh, 0.0, self.dn1, 0.0, g["wg"], g["bg"], "silu", self.space)
        self.dx.copyFrom(c, self.dres)  # the residual's way past the layer; the layer's own share is added to it
        ml.layerNormBackward(c, self.x, p["w1"], self.dn1, 1.0, self.dx, 0.0, g["w1"], g["b1"], self.space, EPSILON)

    def results(self):
        return [self.loss, self.dx] + [self.g[k] for k in sorted(self.g)]


def exact(x, targets, dloss, p):
    n1 = R.layer_norm(x, p["w1"], p["b1"], EPSILON)
    h, kept = R.gated(n1, p["wg"], p["bg"], "silu")
    res = x + h @ p["wd"].T
    n2 = R.layer_norm(res, p["w2"], p["b2"], EPSILON)
    loss = R.cross_entropy(n2, p["wc"], p["bc"], targets)[0]
    g = {}
    dn2, g["wc"], g["bc"] = R.cross_entropy_gradients(n2, p["wc"], p["bc"], targets, dloss)
    dres, g["w2"], g["b2"] = R.layer_norm_gradients(res, p["w2"], dn2, EPSILON)
    g["wd"] = dres.T @ h
    dn1, g["wg"], g["bg"] = R.gated_gradients(n1, p["wg"], kept, dres @ p["wd"], "silu")
    dx, g["w1"], g["b1"] = R.layer_norm_gradients(x, p["w1"], dn1, EPSILON)
    return [loss, dres + dx] + [g[k] for k in sorted(g)]


def case(dtype, rows, features, hidden, classes, seed=1):
    rng = np.random.default_rng(seed)
    p = parameters(rng, features, hidden, classes)
    x, targets = rng.standard_normal((rows, features)), rng.integers(0, classes, rows).astype(np.int32)
    targets[::7] = -1
    dloss = np.full(rows, 0.5, np.float32)
    stored = lambda a: R.numbers(R.bits(a, dtype))
    return x, targets, dloss, p, stored(x), {k: stored(v) for k, v in p.items()}


@pytest.mark.parametrize("dtype,tolerance", [
    # ten roundings to fp16 lie one behind the other (values of 2^-11 / sqrt 3 each, some towards zero in gemm_ex and gemm: 2^-11), none amplified by more than about 2 in norm: 10 * 2 * 2^-11
    ("float16", 10 * 2 * 2.0 ** -11),
    # the same ten operators in fp32, sums of at most 1500 products, errors growing with the root of that: 10 * 2 * 40 * 2^-24
    ("float32", 10 * 2 * 40 * 2.0 ** -24)])
@pytest.mark.parametrize("rows,features,hidden,classes", [(3, 64, 40, 300), (150, 72, 200, 1500), (700, 33, 64, 130)])
def test_a_training_step(ctx, rows, features, hidden, classes, dtype, tolerance):
    x, targets, dloss, p, xs, ps = case(dtype, rows, features, hidden, classes)
    step = Step(ctx, x, targets, dloss, p, dtype)
    step.forward()
    step.backward()
    for got, want in zip(step.results(), exact(xs, targets, dloss.astype(np.float64), ps)):
        off = np.linalg.norm(R.numbers(got.copyToHost(ctx)) - want) / np.linalg.norm(want)
        assert off <= tolerance


def test_a_recorded_step_and_another_one_beside_it(ctx):
    """Forward and backward as one graph on one stream, while a second context makes its own steps eagerly: the eager bits every time."""
    x, targets, dloss, p, _, _ = case("float16", 300, 128, 96, 2000)
    other = ml.Context(0)
    mine, theirs = Step(ctx, x, targets, dloss, p, "float16"), Step(other, x, targets, dloss, p, "float16")

    def both(step):
        step.forward()
        step.backward()

    both(mine)
    eager = [t.copyToHost(ctx) for t in mine.results()]
    with ml.Graph.record(ctx, lambda: both(mine)) as graph:
        for _ in range(3):
            for t in mine.results():
                t.zeroall(ctx)
            graph.launch()
            both(theirs)
            graph.launch()
            ctx.synchronize()
            other.synchronize()
            for step in (mine, theirs):
                assert all(np.array_equal(t.copyToHost(ctx), e) for t, e in zip(step.results(), eager))
    other.destroy()
