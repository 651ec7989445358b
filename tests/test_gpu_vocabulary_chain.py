"""The embedding, the losses over a vocabulary and their gradients as a program uses them together: tokens go in by the embedding, through a normalisation, and come out as the likelihoods of sampled tokens; a
policy loss and a teacher's distillation teach the same weights, whose gradients and the table's are added up; recorded as a graph, beside another stream, with one workspace for all."""
import numpy as np
import pytest

import training_reference as R
import vocabulary_reference as V
from minml_amd import core as ml

pytestmark = pytest.mark.gpu
EPSILON, CLIP, KL_WEIGHT, TEMPERATURE = 1e-5, (0.2, 0.28), float(np.float32(0.05)), 2.0


class Step:
    """Everything a program keeps, and the calls it makes. The output layer has the embedding's table as its weights: three operators add to the gradient of one table, in fp32."""

    def __init__(self, ctx, data, dtype):
        self.ctx, self.data = ctx, data
        dev = lambda a: ml.toDevice(ctx, a)
        for name in ("tokens", "targets", "old", "reference", "advantages", "named", "taught", "dloss", "dteacher"):
            setattr(self, name, dev(data[name]))
        for name in ("table", "w", "b", "bc"):
            setattr(self, name, dev(R.bits(data[name], dtype)))
        sequences, length = data["tokens"].shape
        classes, features = data["table"].shape
        count = data["named"].shape[-1]
        new = lambda *s, d=dtype: ml.Tensor(s, d)
        self.scale, self.classes = float(np.float32(np.sqrt(features))), classes
        self.x, self.n, self.dn, self.dx = (new(sequences, length, features) for _ in range(4))
        self.nll, self.lse, self.lse_t, self.divergence, self.dnll = (new(sequences, length, d="float32") for _ in range(5))
        self.log_p = new(sequences, length, count, d="float32")
        self.loss, self.weights = new(4, d="float32"), new(sequences, d="float32")
        self.dtable, self.dbc, self.dw, self.db = new(classes, features, d="float32"), new(classes, d="float32"), new(features, d="float32"), new(features, d="float32")
        sizes = [ml.linearCrossEntropyGetWorkspaceSize(ctx, self.n, self.table, True), ml.linearDistillationGetWorkspaceSize(ctx, self.n, self.table, count, True),
                 ml.policyLossGetWorkspaceSize(ctx, self.nll), ml.layerNormGetWorkspaceSize(ctx, self.x), ml.embeddingGetWorkspaceSize(ctx, self.tokens, self.dtable)]
        self.space = new(max(sizes), d="uint8")
        self.space.setall(ctx, 0xff)

    def run(self):
        c, s = self.ctx, self.space
        policy = (self.nll, self.old, self.reference, self.advantages, self.targets, self.classes, CLIP, KL_WEIGHT)
        ml.embeddingForward(c, self.tokens, self.table, self.scale, self.x)
        ml.layerNormForward(c, self.x, self.w, self.b, self.n, EPSILON)
        ml.linearCrossEntropyForward(c, self.n, self.table, self.bc, self.targets, self.nll, self.lse, s)
        ml.policyLossForward(c, *policy, "sequences", self.loss, self.weights, s)
        ml.linearDistillationForward(c, self.n, self.table, self.bc, self.named, self.taught, TEMPERATURE, self.divergence, self.lse_t, self.log_p, s)
        ml.policyLossBackward(c, *policy, self.weights, self.dloss, 0.0, self.dnll)
        ml.linearCrossEntropyBackward(c, self.n, self.table, self.bc, self.targets, self.lse, self.dnll, 0.0, self.dn, 0.0, self.dtable, self.dbc, s)
        ml.linearDistillationBackward(c, self.n, self.table, self.bc, self.named, self.taught, TEMPERATURE, self.lse_t, self.log_p, self.dteacher, 1.0, self.dn, 1.0, self.dtable, self.dbc, s)
        ml.layerNormBackward(c, self.x, self.w, self.dn, 0.0, self.dx, 0.0, self.dw, self.db, s, EPSILON)
        ml.embeddingBackward(c, self.tokens, self.dx, self.scale, 1.0, self.dtable, s)

    def results(self):
        return [self.loss, self.divergence, self.dnll, self.dx, self.dtable, self.dbc, self.dw, self.db]


def exact(d, scale):
    rows = lambda a: a.reshape((-1,) + a.shape[2:])
    tokens, targets, named, taught = (rows(d[k]) for k in ("tokens", "targets", "named", "taught"))
    x = V.embedding(tokens, d["table"], scale)
    n = R.layer_norm(x, d["w"], d["b"], EPSILON)
    nll = R.cross_entropy(n, d["table"], d["bc"], targets)[0].reshape(d["tokens"].shape)
    loss, _, dnll = V.policy(nll, d["old"], d["reference"], d["advantages"], d["targets"], len(d["table"]), CLIP, KL_WEIGHT, "sequences")[0]
    dnll = dnll * d["dloss"][0]
    divergence = V.distillation(n, d["table"], d["bc"], named, taught, TEMPERATURE)[0]
    first = R.cross_entropy_gradients(n, d["table"], d["bc"], targets, dnll.reshape(-1))
    second = V.distillation_gradients(n, d["table"], d["bc"], named, taught, TEMPERATURE, rows(d["dteacher"]))
    dn, dtable, dbc = (a + b for a, b in zip(first, second))
    dx, dw, db = R.layer_norm_gradients(x, d["w"], dn, EPSILON)
    dtable = dtable + V.embedding_gradient(tokens, dx, len(dtable), scale)[0]
    return [loss, divergence, dnll.reshape(-1), dx, dtable, dbc, dw, db]


def case(dtype, sequences, length, features, classes, count, seed=1):
    rng = np.random.default_rng(seed)
    shape = (sequences, length)
    table = rng.standard_normal((classes, features)) / np.sqrt(features)
    targets = rng.integers(0, classes, shape)
    targets[:, :length // 4] = -1
    data = dict(tokens=rng.integers(-1, classes, shape).astype(np.int32), targets=targets.astype(np.int32), table=table, w=1 + 0.1 * rng.standard_normal(features), b=0.1 * rng.standard_normal(features),
                bc=0.1 * rng.standard_normal(classes), advantages=rng.standard_normal(sequences).astype(np.float32),
                named=np.argsort(rng.random((sequences, length, classes)), -1)[..., :count].astype(np.int32), taught=rng.standard_normal((sequences, length, count)).astype(np.float32),
                dloss=np.full(1, 64.0, np.float32), dteacher=np.full(shape, 0.02, np.float32))
    stored = {k: R.numbers(R.bits(v, dtype)) if k in ("table", "w", "b", "bc") else v for k, v in data.items()}
    # the sampled tokens' likelihoods a little off what they are now, so that the clip holds some of them and none is near its border
    n = R.layer_norm(V.embedding(data["tokens"].reshape(-1), stored["table"], float(np.float32(np.sqrt(features)))), stored["w"], stored["b"], EPSILON)
    nll = R.cross_entropy(n, stored["table"], stored["bc"], targets.reshape(-1))[0].reshape(shape)
    data["old"] = (nll + rng.choice([-0.5, -0.1, 0.05, 0.12, 0.4], shape)).astype(np.float32)
    data["reference"] = (nll + rng.normal(0, 0.3, shape)).astype(np.float32)
    for k in ("old", "reference"):
        stored[k] = data[k].astype(np.float64)
    return data, stored


@pytest.mark.parametrize("dtype,tolerance", [
    # six roundings to fp16 lie one behind the other (values of 2^-11 / sqrt 3 each), none amplified by more than about 4 in norm, where both losses' gradients partly cancel: 6 * 4 * 2^-11
    ("float16", 6 * 4 * 2.0 ** -11),
    # the same operators in fp32, sums of at most 1500 products, errors growing with the root of that: 6 * 4 * 40 * 2^-24
    ("float32", 6 * 4 * 40 * 2.0 ** -24)])
@pytest.mark.parametrize("sequences,length,features,classes,count", [(1, 5, 64, 300, 7), (6, 40, 72, 1500, 16), (30, 33, 40, 130, 50)])
def test_a_training_step(ctx, sequences, length, features, classes, count, dtype, tolerance):
    data, stored = case(dtype, sequences, length, features, classes, count)
    step = Step(ctx, data, dtype)
    step.run()
    for got, want in zip(step.results(), exact(stored, step.scale)):
        got = R.numbers(got.copyToHost(ctx)).reshape(want.shape)
        assert np.linalg.norm(got - want) <= tolerance * np.linalg.norm(want)


def test_a_recorded_step_and_another_one_beside_it(ctx):
    """All of it as one graph on one stream, while a second context makes its own steps eagerly, each with a workspace of its own: the eager bits every time, also from a workspace that held something else before."""
    data, _ = case("float16", 8, 1100, 64, 2000, 20)
    other = ml.Context(0)
    mine, theirs = Step(ctx, data, "float16"), Step(other, data, "float16")
    mine.run()
    eager = [t.copyToHost(ctx) for t in mine.results()]
    with ml.Graph.record(ctx, mine.run) as graph:
        for _ in range(3):
            for t in mine.results() + [mine.space]:
                t.setall(ctx, 77)
            graph.launch()
            theirs.run()
            graph.launch()
            ctx.synchronize()
            other.synchronize()
            for step in (mine, theirs):
                assert all(np.array_equal(t.copyToHost(ctx), e) for t, e in zip(step.results(), eager))
    other.destroy()


def test_tables_and_batches_of_more_than_2_31_elements(ctx):
    """Offsets that pass 32 bits: the last rows of a table of 2.9e9 elements, looked up and added to; 2.3e9 tokens of the policy loss."""
    classes, features = 70001, 41000
    table = ml.Tensor((classes, features), "float16")
    table.setall(ctx, 1.5)
    tokens = np.array([classes - 1, 0, classes, classes - 1, 52377], np.int32)
    T, y = ml.toDevice(ctx, tokens), ml.Tensor((5, features), "float16")
    ml.embeddingForward(ctx, T, table, 2.0, y)
    got = R.numbers(y.copyToHost(ctx))
    assert (got[[0, 1, 3, 4]] == 3).all() and (got[2] == 0).all()
    ml.embeddingBackward(ctx, T, y, 0.5, 1.0, table, ml.Tensor((ml.embeddingGetWorkspaceSize(ctx, T, table),), "uint8"))
    for row, want in ((0, 3.0), (1, 1.5), (52377, 3.0), (classes - 2, 1.5), (classes - 1, 4.5)):
        assert (R.numbers(table.view((features,), row * features).copyToHost(ctx)) == want).all()
    # every row of dy names the table's last class or none; the rows of dy itself lie beyond 2^31 elements
    rows = 55000
    ids = np.full(rows, -1, np.int32)
    ids[-3:] = 7
    small = ml.Tensor((9, features), "float32")
    T = ml.toDevice(ctx, ids)
    ml.embeddingBackward(ctx, T, table.view((rows, features)), 1.0, 0.0, small, ml.Tensor((ml.embeddingGetWorkspaceSize(ctx, T, small),), "uint8"))
    got = small.copyToHost(ctx)
    assert (got[7] == 4.5).all() and (np.delete(got, 7, 0) == 0).all()
    del table, small, y
    sequences, length = 60001, 38000
    nll, old, dnll = (ml.Tensor((sequences, length), "float32") for _ in range(3))
    targets = ml.Tensor((sequences, length), "int32")
    nll.setall(ctx, 1.0)
    old.setall(ctx, 1.0)
    targets.setall(ctx, -1)
    targets.view((length,), (sequences - 1) * length).setall(ctx, 3)
    loss, weights = ml.Tensor((4,), "float32"), ml.Tensor((sequences,), "float32")
    advantages = ml.Tensor((sequences,), "float32")
    advantages.setall(ctx, 2.0)
    space = ml.Tensor((ml.policyLossGetWorkspaceSize(ctx, nll),), "uint8")
    ml.policyLossForward(ctx, nll, old, None, advantages, targets, 10, (0.2, 0.2), 0.0, "tokens", loss, weights, space)
    assert np.array_equal(loss.copyToHost(ctx), np.array([-2, -2, 0, 0], np.float32))
    assert weights.copyToHost(ctx)[-1] == np.float32(1 / length) and (weights.copyToHost(ctx)[:-1] == 0).all()
    ml.policyLossBackward(ctx, nll, old, None, advantages, targets, 10, (0.2, 0.2), 0.0, weights, None, 0.0, dnll)
    assert (dnll.view((length,), (sequences - 1) * length).copyToHost(ctx) == np.float32(2 * np.float32(1 / length))).all() and (dnll.view((2 * length,), (sequences - 3) * length).copyToHost(ctx) == 0).all()
